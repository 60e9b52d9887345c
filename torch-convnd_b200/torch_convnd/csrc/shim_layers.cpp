// PyTorch dispatcher kernels of the layer operators: torch_convnd::layer_norm, linear and
// gated_recurrence, their training forms (which also return what the backward needs) and
// their backward operators, over the C ABI of convnd_b200_layers.h.
//
// The differentiable entry points register a C++ autograd function: a training step of a
// small layer is bound by host time, of which a Python formula would take most. The CPU
// kernels validate like the CUDA ones and then refuse.
#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "convnd_b200_layers.h"

namespace convnd_b200 {
namespace {

using OptTensor = std::optional<at::Tensor>;
using Grads = std::tuple<OptTensor, OptTensor, OptTensor>;
using Mask = std::array<bool, 3>;

int32_t dtype_code(at::ScalarType type) {
  switch (type) {
    case at::kHalf:
      return CND_F16;
    case at::kBFloat16:
      return CND_BF16;
    case at::kFloat:
      return CND_F32;
    case at::kDouble:
      return CND_F64;
    default:
      return -1;
  }
}

void check_status(int status) { TORCH_CHECK(status == CND_OK, cnd_last_error()); }

void* current_stream(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// The type of row statistics and carried states: float32, float64 for float64.
at::ScalarType wide_type(const at::Tensor& t) {
  return t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
}

at::Tensor workspace_tensor(size_t bytes, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

void* data_or_null(const OptTensor& t) {
  return t.has_value() && t->defined() ? const_cast<void*>(t->const_data_ptr()) : nullptr;
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void check_input(const char* op, const at::Tensor& input) {
  TORCH_CHECK(input.layout() == at::kStrided, op, " requires strided tensors");
  TORCH_CHECK(input.device().is_cpu() || input.device().is_cuda(), op,
              " supports CPU and CUDA tensors");
  TORCH_CHECK(dtype_code(input.scalar_type()) >= 0, op,
              " supports float16, bfloat16, float32 and float64");
}

void check_like(const char* op, const char* name, const at::Tensor& t, const at::Tensor& input) {
  TORCH_CHECK(t.layout() == at::kStrided && t.device() == input.device() &&
                  t.scalar_type() == input.scalar_type(),
              op, ": ", name, " must have the input's device and dtype");
}

// The tensor as rows of its last dimension, unit stride inside a row and one stride between
// rows: itself when its strides allow that, else a contiguous copy.
struct Rows {
  at::Tensor tensor;
  int64_t stride;
};

Rows as_rows(const at::Tensor& t) {
  const int64_t last = t.dim() - 1;
  const int64_t width = t.size(last);
  if (t.is_contiguous() || t.numel() == 0) return {t, width};
  bool regular = t.stride(last) == 1 || width == 1;
  int64_t stride = 0, expected = 0;
  for (int64_t d = last - 1; d >= 0 && regular; --d) {
    if (t.size(d) == 1) continue;
    if (stride == 0) {
      stride = t.stride(d);
      regular = stride >= width;
    } else {
      regular = t.stride(d) == expected;
    }
    expected = t.stride(d) * t.size(d);
  }
  if (!regular) return {t.contiguous(), width};
  return {t, stride == 0 ? width : stride};
}

// A copy where the data does not start on a 16-byte boundary.
at::Tensor aligned(const at::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 ? t : t.clone();
}

int64_t leading(const at::Tensor& t) {
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
  return rows;
}

[[noreturn]] void refuse_cpu(const char* op) {
  TORCH_CHECK(false, "torch_convnd B200 build: ", op,
              " runs on CUDA devices only; move the tensors to a CUDA device");
}

// First-order gradients only: differentiating them again raises instead of silently giving
// zeros.
torch::autograd::variable_list once_differentiable(const char* op,
                                                   torch::autograd::variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads) {
    if (g.defined()) g = g.detach().requires_grad_(true);
  }
  torch::autograd::DelayedError error(
      std::string("torch_convnd::") + op + " has no second derivative", grads.size());
  return error(std::move(grads));
}

// Whether the backward has to fill the gradient of the i-th tensor argument; arguments that
// are absent have no edge.
struct Edges {
  torch::autograd::AutogradContext* ctx;
  size_t next = 0;
  bool operator()(bool present) { return present && ctx->needs_input_grad(next++); }
};

// Whether a backward may follow. A tangent (forward-mode differentiation) would be lost below the
// autograd key without a word, so it is refused.
bool wants_grad(const char* op, std::initializer_list<const at::Tensor*> tensors) {
  bool wanted = false;
  for (const at::Tensor* t : tensors) {
    if (t == nullptr || !t->defined()) continue;
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "torch_convnd::", op,
                                " does not support forward-mode differentiation");
    wanted = wanted || t->requires_grad();
  }
  return wanted && at::GradMode::is_enabled();
}

const at::Tensor* pointer(const OptTensor& t) { return given(t) ? &*t : nullptr; }
at::Tensor tensor(const OptTensor& t) { return given(t) ? *t : at::Tensor(); }
OptTensor optional(const at::Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// ---- layer norm ------------------------------------------------------------------------

void check_norm(const at::Tensor& input, const OptTensor& weight, const OptTensor& bias) {
  check_input("layer_norm", input);
  TORCH_CHECK(input.dim() >= 1 && input.size(-1) > 0,
              "layer_norm requires a last dimension of at least one element");
  at::ScalarType type = input.scalar_type();
  bool seen = false;
  for (const OptTensor* p : {&weight, &bias}) {
    if (!given(*p)) continue;
    TORCH_CHECK((*p)->layout() == at::kStrided && (*p)->dim() == 1 &&
                    (*p)->size(0) == input.size(-1) && (*p)->device() == input.device(),
                "layer_norm: weight and bias must be vectors of the last dimension's size on "
                "the input's device");
    TORCH_CHECK((*p)->scalar_type() == input.scalar_type() ||
                    ((*p)->scalar_type() == at::kFloat && input.scalar_type() != at::kDouble),
                "layer_norm: weight and bias must have the input's dtype or float32");
    TORCH_CHECK(!seen || (*p)->scalar_type() == type,
                "layer_norm: weight and bias must have the same dtype");
    type = (*p)->scalar_type();
    seen = true;
  }
}

int32_t param_code(const at::Tensor& input, const OptTensor& weight, const OptTensor& bias) {
  if (given(weight)) return dtype_code(weight->scalar_type());
  if (given(bias)) return dtype_code(bias->scalar_type());
  return dtype_code(input.scalar_type());
}

std::tuple<at::Tensor, at::Tensor> norm_forward(const at::Tensor& input, const OptTensor& weight,
                                                const OptTensor& bias, double eps, bool train) {
  check_norm(input, weight, bias);
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows x = as_rows(input);
  const int64_t rows = leading(input);
  OptTensor w, b;
  if (given(weight)) w = weight->contiguous();
  if (given(bias)) b = bias->contiguous();
  at::Tensor output = at::empty(input.sizes(), input.options());
  at::Tensor stats = at::empty({train ? 2 : 0, rows}, input.options().dtype(wide_type(input)));
  check_status(cnd_layer_norm_forward(
      dtype_code(input.scalar_type()), param_code(input, weight, bias), rows, input.size(-1),
      x.stride, eps, x.tensor.const_data_ptr(), data_or_null(w), data_or_null(b),
      output.mutable_data_ptr(), train ? stats.mutable_data_ptr() : nullptr,
      current_stream(input)));
  return {output, stats};
}

at::Tensor layer_norm_cuda(const at::Tensor& input, const OptTensor& weight,
                           const OptTensor& bias, double eps) {
  return std::get<0>(norm_forward(input, weight, bias, eps, false));
}

std::tuple<at::Tensor, at::Tensor> layer_norm_train_cuda(const at::Tensor& input,
                                                         const OptTensor& weight,
                                                         const OptTensor& bias, double eps) {
  return norm_forward(input, weight, bias, eps, true);
}

void check_norm_backward(const at::Tensor& grad_output, const at::Tensor& input,
                         const OptTensor& weight, const OptTensor& bias,
                         const at::Tensor& stats) {
  check_norm(input, weight, bias);
  check_like("layer_norm_backward", "grad_output", grad_output, input);
  TORCH_CHECK(grad_output.sizes() == input.sizes(),
              "layer_norm_backward: grad_output must have the input's shape");
  TORCH_CHECK(stats.layout() == at::kStrided && stats.device() == input.device() &&
                  stats.scalar_type() == wide_type(input) && stats.is_contiguous() &&
                  stats.dim() == 2 && stats.size(0) == 2 && stats.size(1) == leading(input),
              "layer_norm_backward: stats must be the statistics of the input's rows");
}

Grads layer_norm_backward_cuda(const at::Tensor& grad_output, const at::Tensor& input,
                               const OptTensor& weight, const OptTensor& bias,
                               const at::Tensor& stats, Mask output_mask) {
  check_norm_backward(grad_output, input, weight, bias, stats);
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows x = as_rows(input), dy = as_rows(grad_output);
  const int64_t rows = leading(input), width = input.size(-1);
  OptTensor w, dx, dweight, dbias;
  if (given(weight)) w = weight->contiguous();
  const at::TensorOptions params =
      input.options().dtype(given(weight) ? weight->scalar_type()
                                          : given(bias) ? bias->scalar_type()
                                                        : input.scalar_type());
  if (output_mask[0]) dx = at::empty(input.sizes(), input.options());
  if (output_mask[1]) dweight = at::empty({width}, params);
  if (output_mask[2]) dbias = at::empty({width}, params);
  const int32_t mask[3] = {output_mask[0], output_mask[1], output_mask[2]};
  const int32_t dtype = dtype_code(input.scalar_type());
  const size_t bytes = cnd_layer_norm_backward_workspace_size(dtype, rows, width, mask);
  at::Tensor workspace = workspace_tensor(bytes, input);
  check_status(cnd_layer_norm_backward(
      dtype, param_code(input, weight, bias), rows, width, dy.stride, x.stride,
      dy.tensor.const_data_ptr(), x.tensor.const_data_ptr(), data_or_null(w),
      stats.const_data_ptr(), data_or_null(dx), data_or_null(dweight), data_or_null(dbias), mask,
      workspace.mutable_data_ptr(), bytes, current_stream(input)));
  return {dx, dweight, dbias};
}

at::Tensor layer_norm_cpu(const at::Tensor& input, const OptTensor& weight, const OptTensor& bias,
                          double eps) {
  (void)eps;
  check_norm(input, weight, bias);
  refuse_cpu("layer_norm");
}

std::tuple<at::Tensor, at::Tensor> layer_norm_train_cpu(const at::Tensor& input,
                                                        const OptTensor& weight,
                                                        const OptTensor& bias, double eps) {
  (void)eps;
  check_norm(input, weight, bias);
  refuse_cpu("layer_norm");
}

Grads layer_norm_backward_cpu(const at::Tensor& grad_output, const at::Tensor& input,
                              const OptTensor& weight, const OptTensor& bias,
                              const at::Tensor& stats, Mask output_mask) {
  (void)output_mask;
  check_norm_backward(grad_output, input, weight, bias, stats);
  refuse_cpu("layer_norm");
}

template <typename Signature>
c10::TypedOperatorHandle<Signature> find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

class LayerNormFunction : public torch::autograd::Function<LayerNormFunction> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& input,
                            const OptTensor& weight, const OptTensor& bias, double eps) {
    static const auto op =
        find_op<decltype(layer_norm_train_cuda)>("torch_convnd::layer_norm_train");
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [output, stats] = op.call(input, weight, bias, eps);
    ctx->save_for_backward({input, tensor(weight), tensor(bias), stats});
    return output;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    static const auto op =
        find_op<decltype(layer_norm_backward_cuda)>("torch_convnd::layer_norm_backward");
    const auto saved = ctx->get_saved_variables();
    Edges needs{ctx};
    const bool dx = needs(true), dw = needs(saved[1].defined()), db = needs(saved[2].defined());
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto [gx, gw, gb] = op.call(grads[0], saved[0], optional(saved[1]), optional(saved[2]),
                                      saved[3], Mask{dx, dw, db});
    return once_differentiable("layer_norm", {tensor(gx), tensor(gw), tensor(gb), at::Tensor()});
  }
};

at::Tensor layer_norm_autograd(const at::Tensor& input, const OptTensor& weight,
                               const OptTensor& bias, double eps) {
  if (wants_grad("layer_norm", {&input, pointer(weight), pointer(bias)})) {
    return LayerNormFunction::apply(input, weight, bias, eps);
  }
  static const auto op = find_op<decltype(layer_norm_cuda)>("torch_convnd::layer_norm");
  at::AutoDispatchBelowADInplaceOrView guard;
  return op.call(input, weight, bias, eps);
}

// ---- linear ----------------------------------------------------------------------------

int32_t activation_code(c10::string_view activation) {
  if (activation == "none") return CND_ACT_NONE;
  if (activation == "gelu") return CND_ACT_GELU;
  if (activation == "silu") return CND_ACT_SILU;
  TORCH_CHECK(false, "linear supports activation='none', 'gelu' or 'silu', got '",
              std::string(activation), "'");
}

std::vector<int64_t> linear_shape(const at::Tensor& input, const at::Tensor& weight) {
  std::vector<int64_t> shape = input.sizes().vec();
  shape.back() = weight.size(0);
  return shape;
}

cnd_linear check_linear(const at::Tensor& input, const at::Tensor& weight, const OptTensor& bias,
                        const OptTensor& residual, c10::string_view activation) {
  cnd_linear p{};
  p.activation = activation_code(activation);
  check_input("linear", input);
  check_like("linear", "weight", weight, input);
  TORCH_CHECK(input.dim() >= 1 && weight.dim() == 2 && weight.size(1) == input.size(-1) &&
                  weight.size(0) > 0 && weight.size(1) > 0,
              "linear: weight must be [out_features, in_features] with the input's last "
              "dimension as in_features, both positive");
  if (given(bias)) {
    check_like("linear", "bias", *bias, input);
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0),
                "linear: bias must be a vector of out_features");
  }
  if (given(residual)) {
    check_like("linear", "residual", *residual, input);
    TORCH_CHECK(residual->sizes() == at::IntArrayRef(linear_shape(input, weight)),
                "linear: residual must have the output's shape");
  }
  p.dtype = dtype_code(input.scalar_type());
  p.rows = leading(input);
  p.in_features = weight.size(1);
  p.out_features = weight.size(0);
  p.x_stride = p.in_features;
  return p;
}

std::tuple<at::Tensor, at::Tensor> linear_forward(const at::Tensor& input,
                                                  const at::Tensor& weight, const OptTensor& bias,
                                                  const OptTensor& residual,
                                                  c10::string_view activation, bool train) {
  cnd_linear p = check_linear(input, weight, bias, residual, activation);
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows x = as_rows(aligned(input));
  p.x_stride = x.stride;
  const at::Tensor w = aligned(weight.contiguous());
  OptTensor b, r;
  if (given(bias)) b = bias->contiguous();
  if (given(residual)) r = residual->contiguous();
  const std::vector<int64_t> shape = linear_shape(input, weight);
  at::Tensor output = at::empty(shape, input.options());
  const bool keep = train && p.activation != CND_ACT_NONE;
  at::Tensor pre = keep ? at::empty(shape, input.options()) : at::empty({0}, input.options());
  const size_t bytes = cnd_linear_forward_workspace_size(&p);
  at::Tensor workspace;
  if (bytes > 0) workspace = workspace_tensor(bytes, input);
  check_status(cnd_linear_forward(
      &p, x.tensor.const_data_ptr(), w.const_data_ptr(), data_or_null(b), data_or_null(r),
      output.mutable_data_ptr(), keep ? pre.mutable_data_ptr() : nullptr,
      bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, current_stream(input)));
  return {output, pre};
}

at::Tensor linear_cuda(const at::Tensor& input, const at::Tensor& weight, const OptTensor& bias,
                       const OptTensor& residual, c10::string_view activation) {
  return std::get<0>(linear_forward(input, weight, bias, residual, activation, false));
}

std::tuple<at::Tensor, at::Tensor> linear_train_cuda(const at::Tensor& input,
                                                     const at::Tensor& weight,
                                                     const OptTensor& bias,
                                                     const OptTensor& residual,
                                                     c10::string_view activation) {
  return linear_forward(input, weight, bias, residual, activation, true);
}

cnd_linear check_linear_backward(const at::Tensor& grad_output, const at::Tensor& pre,
                                 const at::Tensor& input, const at::Tensor& weight,
                                 c10::string_view activation) {
  const cnd_linear p = check_linear(input, weight, std::nullopt, std::nullopt, activation);
  const std::vector<int64_t> shape = linear_shape(input, weight);
  check_like("linear_backward", "grad_output", grad_output, input);
  check_like("linear_backward", "pre", pre, input);
  TORCH_CHECK(grad_output.sizes() == at::IntArrayRef(shape),
              "linear_backward: grad_output must have the output's shape");
  TORCH_CHECK(p.activation == CND_ACT_NONE || pre.sizes() == at::IntArrayRef(shape),
              "linear_backward: pre must have the output's shape");
  return p;
}

Grads linear_backward_cuda(const at::Tensor& grad_output, const at::Tensor& pre,
                           const at::Tensor& input, const at::Tensor& weight,
                           c10::string_view activation, Mask output_mask) {
  cnd_linear p = check_linear_backward(grad_output, pre, input, weight, activation);
  const c10::cuda::CUDAGuard guard(input.device());
  const Rows x = as_rows(aligned(input));
  p.x_stride = x.stride;
  const at::Tensor dy = aligned(grad_output.contiguous()), w = aligned(weight.contiguous());
  const at::Tensor z = aligned(pre.contiguous());
  OptTensor dx, dweight, dbias;
  if (output_mask[0]) dx = at::empty(input.sizes(), input.options());
  if (output_mask[1]) dweight = at::empty(weight.sizes(), weight.options());
  if (output_mask[2]) dbias = at::empty({weight.size(0)}, weight.options());
  const int32_t mask[3] = {output_mask[0], output_mask[1], output_mask[2]};
  const size_t bytes = cnd_linear_backward_workspace_size(&p, mask);
  at::Tensor workspace;
  if (bytes > 0) workspace = workspace_tensor(bytes, input);
  check_status(cnd_linear_backward(
      &p, dy.const_data_ptr(), p.activation == CND_ACT_NONE ? nullptr : z.const_data_ptr(),
      x.tensor.const_data_ptr(), w.const_data_ptr(), data_or_null(dx), data_or_null(dweight),
      data_or_null(dbias), mask, bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes,
      current_stream(input)));
  return {dx, dweight, dbias};
}

at::Tensor linear_cpu(const at::Tensor& input, const at::Tensor& weight, const OptTensor& bias,
                      const OptTensor& residual, c10::string_view activation) {
  check_linear(input, weight, bias, residual, activation);
  refuse_cpu("linear");
}

std::tuple<at::Tensor, at::Tensor> linear_train_cpu(const at::Tensor& input,
                                                    const at::Tensor& weight,
                                                    const OptTensor& bias,
                                                    const OptTensor& residual,
                                                    c10::string_view activation) {
  check_linear(input, weight, bias, residual, activation);
  refuse_cpu("linear");
}

Grads linear_backward_cpu(const at::Tensor& grad_output, const at::Tensor& pre,
                          const at::Tensor& input, const at::Tensor& weight,
                          c10::string_view activation, Mask output_mask) {
  (void)output_mask;
  check_linear_backward(grad_output, pre, input, weight, activation);
  refuse_cpu("linear");
}

class LinearFunction : public torch::autograd::Function<LinearFunction> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& input,
                            const at::Tensor& weight, const OptTensor& bias,
                            const OptTensor& residual, c10::string_view activation) {
    static const auto op = find_op<decltype(linear_train_cuda)>("torch_convnd::linear_train");
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [output, pre] = op.call(input, weight, bias, residual, activation);
    ctx->save_for_backward({input, weight, pre});
    ctx->saved_data["activation"] = std::string(activation);
    ctx->saved_data["bias"] = given(bias);
    ctx->saved_data["residual"] = given(residual);
    return output;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    static const auto op =
        find_op<decltype(linear_backward_cuda)>("torch_convnd::linear_backward");
    const auto saved = ctx->get_saved_variables();
    Edges needs{ctx};
    const bool dx = needs(true), dw = needs(true);
    const bool db = needs(ctx->saved_data["bias"].toBool());
    const bool dr = needs(ctx->saved_data["residual"].toBool());
    at::AutoDispatchBelowADInplaceOrView guard;
    Grads g;
    if (dx || dw || db) {
      g = op.call(grads[0], saved[2], saved[0], saved[1],
                  ctx->saved_data["activation"].toStringRef(), Mask{dx, dw, db});
    }
    return once_differentiable(
        "linear", {tensor(std::get<0>(g)), tensor(std::get<1>(g)), tensor(std::get<2>(g)),
                   dr ? grads[0] : at::Tensor(), at::Tensor()});
  }
};

at::Tensor linear_autograd(const at::Tensor& input, const at::Tensor& weight,
                           const OptTensor& bias, const OptTensor& residual,
                           c10::string_view activation) {
  if (wants_grad("linear", {&input, &weight, pointer(bias), pointer(residual)})) {
    return LinearFunction::apply(input, weight, bias, residual, activation);
  }
  static const auto op = find_op<decltype(linear_cuda)>("torch_convnd::linear");
  at::AutoDispatchBelowADInplaceOrView guard;
  return op.call(input, weight, bias, residual, activation);
}

template <c10::DeviceType Device>
at::Tensor linear_autocast(const at::Tensor& input, const at::Tensor& weight,
                           const OptTensor& bias, const OptTensor& residual,
                           c10::string_view activation) {
  const c10::impl::ExcludeDispatchKeyGuard no_autocast(
      at::autocast::get_autocast_dispatch_key_from_device_type(Device));
  const at::ScalarType target = at::autocast::get_autocast_dtype(Device);
  static const auto op = find_op<decltype(linear_cuda)>("torch_convnd::linear");
  return op.call(at::autocast::cached_cast(target, input, Device),
                 at::autocast::cached_cast(target, weight, Device),
                 at::autocast::cached_cast(target, bias, Device),
                 at::autocast::cached_cast(target, residual, Device), activation);
}

// ---- gated recurrence ------------------------------------------------------------------

// A dense tensor in memory order: `outer` x `steps` x `inner` around the recurrence's axis,
// and the sizes and strides of a state (the tensor without that axis, same memory order).
struct Columns {
  at::Tensor x;
  int64_t outer = 1, steps = 0, inner = 1;
  std::vector<int64_t> state_sizes, state_strides;
};

int64_t check_recurrence(const at::Tensor& input, const at::Tensor& gate, const OptTensor& initial,
                         int64_t dim) {
  check_input("gated_recurrence", input);
  TORCH_CHECK(input.dim() >= 1 && dim >= -input.dim() && dim < input.dim(),
              "gated_recurrence: dim must be a dimension of the input");
  dim = dim < 0 ? dim + input.dim() : dim;
  check_like("gated_recurrence", "gate", gate, input);
  TORCH_CHECK(gate.sizes() == input.sizes(), "gated_recurrence: gate must have the input's shape");
  if (given(initial)) {
    std::vector<int64_t> state = input.sizes().vec();
    state.erase(state.begin() + dim);
    TORCH_CHECK(initial->layout() == at::kStrided && initial->device() == input.device() &&
                    initial->scalar_type() == wide_type(input) &&
                    initial->sizes() == at::IntArrayRef(state),
                "gated_recurrence: initial must be the input's shape without dim, float32 "
                "(float64 for a float64 input), on the input's device");
  }
  return dim;
}

Columns columns_of(const at::Tensor& input, int64_t dim) {
  Columns c;
  c.x = input.is_non_overlapping_and_dense() ? input : input.contiguous();
  c.steps = input.size(dim);
  const int64_t own = c.x.stride(dim);
  for (int64_t d = 0; d < input.dim(); ++d) {
    if (d == dim) continue;
    const int64_t size = input.size(d), stride = c.x.stride(d);
    // with at most one step no axis lies outside it
    const bool outside = c.steps > 1 && size > 1 && stride > own;
    (outside ? c.outer : c.inner) *= size;
    c.state_sizes.push_back(size);
    c.state_strides.push_back(outside ? stride / c.steps : stride);
  }
  if (input.numel() == 0) {
    // an empty tensor counts as dense whatever its strides (a slice without steps keeps its
    // source's), so they say nothing about a dense state
    int64_t next = 1;
    for (size_t d = c.state_sizes.size(); d-- > 0;) {
      c.state_strides[d] = next;
      next *= std::max<int64_t>(c.state_sizes[d], 1);
    }
  }
  return c;
}

bool same_strides(const at::Tensor& t, at::IntArrayRef strides) {
  for (int64_t d = 0; d < t.dim(); ++d) {
    if (t.size(d) != 1 && t.stride(d) != strides[d]) return false;
  }
  return true;
}

// `t` with the given strides: itself, or a copy.
at::Tensor with_strides(const at::Tensor& t, at::IntArrayRef strides) {
  if (same_strides(t, strides)) return t;
  at::Tensor copy = at::empty_strided(t.sizes(), strides, t.options());
  copy.copy_(t);
  return copy;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> recurrence_forward(
    const at::Tensor& input, const at::Tensor& gate, const OptTensor& initial, int64_t dim,
    bool train) {
  dim = check_recurrence(input, gate, initial, dim);
  const c10::cuda::CUDAGuard guard(input.device());
  const Columns c = columns_of(input, dim);
  const at::Tensor g = with_strides(gate, c.x.strides());
  OptTensor h0;
  if (given(initial)) h0 = with_strides(*initial, c.state_strides);
  const at::TensorOptions wide = input.options().dtype(wide_type(input));
  at::Tensor output = at::empty_strided(input.sizes(), c.x.strides(), input.options());
  at::Tensor last = at::empty_strided(c.state_sizes, c.state_strides, wide);
  const int32_t dtype = dtype_code(input.scalar_type());
  const int64_t blocks =
      train ? cnd_gated_recurrence_blocks(dtype, c.outer, c.steps, c.inner) : 0;
  at::Tensor states = at::empty({blocks, c.outer * c.inner}, wide);
  const size_t bytes = cnd_gated_recurrence_workspace_size(dtype, c.outer, c.steps, c.inner);
  at::Tensor workspace;
  if (bytes > 0) workspace = workspace_tensor(bytes, input);
  check_status(cnd_gated_recurrence_forward(
      dtype, c.outer, c.steps, c.inner, c.x.const_data_ptr(), g.const_data_ptr(),
      data_or_null(h0), output.mutable_data_ptr(), last.mutable_data_ptr(),
      train ? states.mutable_data_ptr() : nullptr,
      bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, current_stream(input)));
  return {output, last, states};
}

std::tuple<at::Tensor, at::Tensor> gated_recurrence_cuda(const at::Tensor& input,
                                                         const at::Tensor& gate,
                                                         const OptTensor& initial, int64_t dim) {
  auto [output, last, states] = recurrence_forward(input, gate, initial, dim, false);
  return {output, last};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> gated_recurrence_train_cuda(
    const at::Tensor& input, const at::Tensor& gate, const OptTensor& initial, int64_t dim) {
  return recurrence_forward(input, gate, initial, dim, true);
}

int64_t check_recurrence_backward(const OptTensor& grad_output, const OptTensor& grad_last,
                                  const at::Tensor& input, const at::Tensor& gate,
                                  const at::Tensor& states, int64_t dim) {
  dim = check_recurrence(input, gate, grad_last, dim);
  if (given(grad_output)) {
    check_like("gated_recurrence_backward", "grad_output", *grad_output, input);
    TORCH_CHECK(grad_output->sizes() == input.sizes(),
                "gated_recurrence_backward: grad_output must have the input's shape");
  }
  TORCH_CHECK(states.layout() == at::kStrided && states.device() == input.device() &&
                  states.scalar_type() == wide_type(input) && states.is_contiguous() &&
                  states.dim() == 2,
              "gated_recurrence_backward: states must be the forward's states");
  return dim;
}

Grads gated_recurrence_backward_cuda(const OptTensor& grad_output, const OptTensor& grad_last,
                                     const at::Tensor& input, const at::Tensor& gate,
                                     const at::Tensor& states, int64_t dim, Mask output_mask) {
  dim = check_recurrence_backward(grad_output, grad_last, input, gate, states, dim);
  const c10::cuda::CUDAGuard guard(input.device());
  const Columns c = columns_of(input, dim);
  const int32_t dtype = dtype_code(input.scalar_type());
  TORCH_CHECK(states.size(0) == cnd_gated_recurrence_blocks(dtype, c.outer, c.steps, c.inner) &&
                  states.size(1) == c.outer * c.inner,
              "gated_recurrence_backward: states must be the forward's states");
  const at::Tensor g = with_strides(gate, c.x.strides());
  OptTensor dy, dlast, dx, dgate, dinitial;
  if (given(grad_output)) dy = with_strides(*grad_output, c.x.strides());
  if (given(grad_last)) dlast = with_strides(*grad_last, c.state_strides);
  if (output_mask[0]) dx = at::empty_strided(input.sizes(), c.x.strides(), input.options());
  if (output_mask[1]) dgate = at::empty_strided(input.sizes(), c.x.strides(), input.options());
  if (output_mask[2]) {
    dinitial = at::empty_strided(c.state_sizes, c.state_strides,
                                 input.options().dtype(wide_type(input)));
  }
  const int32_t mask[3] = {output_mask[0], output_mask[1], output_mask[2]};
  const size_t bytes = cnd_gated_recurrence_workspace_size(dtype, c.outer, c.steps, c.inner);
  at::Tensor workspace;
  if (bytes > 0) workspace = workspace_tensor(bytes, input);
  check_status(cnd_gated_recurrence_backward(
      dtype, c.outer, c.steps, c.inner, data_or_null(dy), data_or_null(dlast),
      c.x.const_data_ptr(), g.const_data_ptr(), states.const_data_ptr(), data_or_null(dx),
      data_or_null(dgate), data_or_null(dinitial), mask,
      bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, current_stream(input)));
  return {dx, dgate, dinitial};
}

std::tuple<at::Tensor, at::Tensor> gated_recurrence_cpu(const at::Tensor& input,
                                                        const at::Tensor& gate,
                                                        const OptTensor& initial, int64_t dim) {
  check_recurrence(input, gate, initial, dim);
  refuse_cpu("gated_recurrence");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> gated_recurrence_train_cpu(
    const at::Tensor& input, const at::Tensor& gate, const OptTensor& initial, int64_t dim) {
  check_recurrence(input, gate, initial, dim);
  refuse_cpu("gated_recurrence");
}

Grads gated_recurrence_backward_cpu(const OptTensor& grad_output, const OptTensor& grad_last,
                                    const at::Tensor& input, const at::Tensor& gate,
                                    const at::Tensor& states, int64_t dim, Mask output_mask) {
  (void)output_mask;
  check_recurrence_backward(grad_output, grad_last, input, gate, states, dim);
  refuse_cpu("gated_recurrence");
}

class RecurrenceFunction : public torch::autograd::Function<RecurrenceFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const at::Tensor& input, const at::Tensor& gate,
                                                const OptTensor& initial, int64_t dim) {
    static const auto op =
        find_op<decltype(gated_recurrence_train_cuda)>("torch_convnd::gated_recurrence_train");
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [output, last, states] = op.call(input, gate, initial, dim);
    ctx->save_for_backward({input, gate, states});
    ctx->saved_data["dim"] = dim;
    ctx->saved_data["initial"] = given(initial);
    // an output that the loss does not use sends no gradient, not a tensor of zeros
    ctx->set_materialize_grads(false);
    return {output, last};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    static const auto op = find_op<decltype(gated_recurrence_backward_cuda)>(
        "torch_convnd::gated_recurrence_backward");
    const auto saved = ctx->get_saved_variables();
    Edges needs{ctx};
    const bool dx = needs(true), dg = needs(true);
    const bool d0 = needs(ctx->saved_data["initial"].toBool());
    if (!grads[0].defined() && !grads[1].defined()) return {{}, {}, {}, {}};
    at::AutoDispatchBelowADInplaceOrView guard;
    const auto [gx, gg, g0] =
        op.call(optional(grads[0]), optional(grads[1]), saved[0], saved[1], saved[2],
                ctx->saved_data["dim"].toInt(), Mask{dx, dg, d0});
    return once_differentiable("gated_recurrence",
                               {tensor(gx), tensor(gg), tensor(g0), at::Tensor()});
  }
};

std::tuple<at::Tensor, at::Tensor> gated_recurrence_autograd(const at::Tensor& input,
                                                             const at::Tensor& gate,
                                                             const OptTensor& initial,
                                                             int64_t dim) {
  if (wants_grad("gated_recurrence", {&input, &gate, pointer(initial)})) {
    auto outputs = RecurrenceFunction::apply(input, gate, initial, dim);
    return {outputs[0], outputs[1]};
  }
  static const auto op = find_op<decltype(gated_recurrence_cuda)>("torch_convnd::gated_recurrence");
  at::AutoDispatchBelowADInplaceOrView guard;
  return op.call(input, gate, initial, dim);
}

}  // namespace
}  // namespace convnd_b200

TORCH_LIBRARY_IMPL(torch_convnd, CUDA, library) {
  library.impl("layer_norm", &convnd_b200::layer_norm_cuda);
  library.impl("layer_norm_train", &convnd_b200::layer_norm_train_cuda);
  library.impl("layer_norm_backward", &convnd_b200::layer_norm_backward_cuda);
  library.impl("linear", &convnd_b200::linear_cuda);
  library.impl("linear_train", &convnd_b200::linear_train_cuda);
  library.impl("linear_backward", &convnd_b200::linear_backward_cuda);
  library.impl("gated_recurrence", &convnd_b200::gated_recurrence_cuda);
  library.impl("gated_recurrence_train", &convnd_b200::gated_recurrence_train_cuda);
  library.impl("gated_recurrence_backward", &convnd_b200::gated_recurrence_backward_cuda);
}

TORCH_LIBRARY_IMPL(torch_convnd, CPU, library) {
  library.impl("layer_norm", &convnd_b200::layer_norm_cpu);
  library.impl("layer_norm_train", &convnd_b200::layer_norm_train_cpu);
  library.impl("layer_norm_backward", &convnd_b200::layer_norm_backward_cpu);
  library.impl("linear", &convnd_b200::linear_cpu);
  library.impl("linear_train", &convnd_b200::linear_train_cpu);
  library.impl("linear_backward", &convnd_b200::linear_backward_cpu);
  library.impl("gated_recurrence", &convnd_b200::gated_recurrence_cpu);
  library.impl("gated_recurrence_train", &convnd_b200::gated_recurrence_train_cpu);
  library.impl("gated_recurrence_backward", &convnd_b200::gated_recurrence_backward_cpu);
}

TORCH_LIBRARY_IMPL(torch_convnd, Autograd, library) {
  library.impl("layer_norm", &convnd_b200::layer_norm_autograd);
  library.impl("linear", &convnd_b200::linear_autograd);
  library.impl("gated_recurrence", &convnd_b200::gated_recurrence_autograd);
}

TORCH_LIBRARY_IMPL(torch_convnd, AutocastCUDA, library) {
  library.impl("linear", &convnd_b200::linear_autocast<c10::DeviceType::CUDA>);
}

TORCH_LIBRARY_IMPL(torch_convnd, AutocastCPU, library) {
  library.impl("linear", &convnd_b200::linear_autocast<c10::DeviceType::CPU>);
}
