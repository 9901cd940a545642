// linear: checks, allocation and autograd around rfm_linear_*.
#include <ATen/autocast_mode.h>

#include "host_common.h"

namespace rfm_host {
namespace {

int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }

bool tma_rows(const Tensor& y) {
  return reinterpret_cast<uintptr_t>(y.data_ptr()) % 16 == 0 && (y.size(0) <= 1 || y.stride(0) % 8 == 0);
}

// `x` as a matrix that TMA can read: rows of adjacent elements, 16-byte aligned,
// their stride a multiple of 8 elements.  A view where the layout allows, else a
// copy with padded rows.
Tensor operand(const Tensor& x) {
  const Tensor y = rows_of(x);
  if (y.numel() == 0 || tma_rows(y)) return y;
  const Tensor copy = at::empty({y.size(0), pad8(y.size(1))}, y.options()).narrow(1, 0, y.size(1));
  copy.copy_(y);
  return copy;
}

int64_t operand_stride(const Tensor& y) { return y.size(0) > 1 ? y.stride(0) : pad8(y.size(1)); }

struct Outputs {
  Tensor out, pre;
  Tensor x, weight;  // as the product read them
};

Outputs forward_rows(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t activation,
                     const Tensor& residual, bool keep_pre) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = weight.size(0);
  Outputs o;
  o.out = at::empty(shape, x.options().memory_format(at::MemoryFormat::Contiguous));
  const Tensor xs = operand(x), ws = operand(weight);
  const int64_t rows = xs.size(0);
  o.x = xs;
  o.weight = ws;
  if (keep_pre) o.pre = at::empty({rows, weight.size(0)}, x.options().memory_format(at::MemoryFormat::Contiguous));
  if (rows == 0) return o;
  const Tensor res = residual.defined() ? rows_of(residual) : Tensor();
  rfm_linear a{};
  a.x = xs.data_ptr();
  a.weight = ws.data_ptr();
  a.bias = data_or_null(bias);
  a.residual = data_or_null(res);
  a.out = o.out.data_ptr();
  a.pre = data_or_null(o.pre);
  a.rows = rows;
  a.ld_x = operand_stride(xs);
  a.ld_weight = operand_stride(ws);
  a.ld_residual = res.defined() ? row_stride(res) : 0;
  a.in_features = static_cast<int32_t>(weight.size(1));
  a.out_features = static_cast<int32_t>(weight.size(0));
  a.dtype = dtype_code(x.scalar_type());
  a.bias_dtype = bias.defined() ? dtype_code(bias.scalar_type()) : a.dtype;
  a.activation = static_cast<int32_t>(activation);
  const int64_t size = rfm_linear_forward_workspace_bytes(rows, a.in_features, a.out_features);
  Tensor work;
  if (size > 0) {
    work = at::empty({size}, x.options().dtype(at::kByte));
    a.workspace = work.data_ptr();
    a.workspace_bytes = size;
  }
  check_call("rfm_linear_forward", rfm_linear_forward(&a, current_stream(x.device())));
  return o;
}

struct Linear : torch::autograd::Function<Linear> {
  // what the backward knows about the call beside the saved tensors
  enum { kActivation, kInFeatures, kType, kBiasType, kBias, kResidual, kCallSize };

  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const MaybeTensor& maybe_bias,
                        int64_t activation, const MaybeTensor& maybe_residual) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const Tensor bias = or_undefined(maybe_bias), residual = or_undefined(maybe_residual);
    // what the wanted gradients read, and nothing else: x for the weight's, the weight for x's, the
    // pre-activation for any that passes the activation.  relu's gradient only asks for its sign, which the
    // output has where nothing was added to it
    const bool for_x = x.requires_grad(), for_w = weight.requires_grad();
    const bool acts =
        activation != RFM_ACT_NONE && (for_x || for_w || (bias.defined() && bias.requires_grad()));
    const bool from_out = activation == RFM_ACT_RELU && !residual.defined();
    const Outputs o = forward_rows(x, weight, bias, activation, residual, acts && !from_out);
    variable_list kept{for_w ? x : Tensor(), for_x ? weight : Tensor(),
                       !acts ? Tensor() : from_out ? o.out : o.pre};
    // operands that had to be copied are kept for the backward, beside the tensors that it checks for changes
    const Tensor x_copy = for_w && !o.x.is_alias_of(x) ? o.x : Tensor();
    const Tensor weight_copy = for_x && !o.weight.is_alias_of(weight) ? o.weight : Tensor();
    if (x_copy.defined() || weight_copy.defined()) {
      kept.push_back(x_copy);
      kept.push_back(weight_copy);
    }
    ctx->save_for_backward(std::move(kept));
    std::vector<int64_t> call(kCallSize);
    call[kActivation] = activation;
    call[kInFeatures] = weight.size(1);
    call[kType] = static_cast<int64_t>(x.scalar_type());
    call[kBiasType] = static_cast<int64_t>(bias.defined() ? bias.scalar_type() : x.scalar_type());
    // places among the tensors given (-1: not given), which number the gradients asked for
    call[kBias] = bias.defined() ? 2 : -1;
    call[kResidual] = residual.defined() ? (bias.defined() ? 3 : 2) : -1;
    ctx->saved_data["call"] = std::move(call);
    return o.out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list result(5);
    if (!grads[0].defined()) return result;
    refuse_tangents("linear's gradient", {&grads[0]});
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> call = ctx->saved_data["call"].toIntVector();
    // saved-tensor hooks may have given everything other strides
    const Tensor kept = saved[2].defined() ? saved[2].contiguous() : Tensor();
    const c10::cuda::CUDAGuard guard(grads[0].device());
    {
      at::AutoGradMode off(false);
      const bool need_bias = call[kBias] > 0 && ctx->needs_input_grad(call[kBias]);
      const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
      const int64_t at_res = call[kResidual], in = call[kInFeatures], out = grads[0].size(-1);
      const auto type = static_cast<at::ScalarType>(call[kType]);
      const Tensor dy = grads[0].scalar_type() == type ? grads[0] : grads[0].to(type);
      if (at_res > 0 && ctx->needs_input_grad(at_res)) result[4] = dy;
      if (need_x || need_w || need_bias) {
        const Tensor g = rows_of(dy);
        const bool copies = saved.size() > 3;
        const Tensor xs = !need_w ? Tensor() : operand(copies && saved[3].defined() ? saved[3] : saved[0]);
        const Tensor ws = !need_x ? Tensor() : operand(copies && saved[4].defined() ? saved[4] : saved[1]);
        const auto options = dy.options().memory_format(at::MemoryFormat::Contiguous);
        rfm_linear_grad a{};
        a.rows = g.size(0);
        a.in_features = static_cast<int32_t>(in);
        a.out_features = static_cast<int32_t>(out);
        a.dtype = dtype_code(type);
        a.activation = static_cast<int32_t>(call[kActivation]);
        const auto bias_type = static_cast<at::ScalarType>(call[kBiasType]);
        a.bias_dtype = dtype_code(bias_type);
        if (need_x) {
          std::vector<int64_t> shape = dy.sizes().vec();
          shape.back() = in;
          result[0] = at::empty(shape, options);
        }
        if (need_w) result[1] = at::empty({out, in}, options);
        if (need_bias) result[2] = at::empty({out}, options.dtype(bias_type));
        a.x = data_or_null(xs);
        a.weight = data_or_null(ws);
        a.saved = data_or_null(kept);
        a.grad_out = g.data_ptr();
        a.ld_x = need_w ? operand_stride(xs) : 0;
        a.ld_weight = need_x ? operand_stride(ws) : 0;
        a.ld_grad = operand_stride(g);
        a.grad_x = data_or_null(result[0]);
        a.grad_weight = data_or_null(result[1]);
        a.grad_bias = data_or_null(result[2]);
        Tensor dp, work;
        if ((need_x || need_w) && a.rows > 0 && (a.activation != RFM_ACT_NONE || !tma_rows(g))) {
          a.ld_grad_pre = pad8(out);
          dp = at::empty({a.rows, a.ld_grad_pre}, options);
          a.grad_pre = dp.data_ptr();
        }
        const int64_t size = rfm_linear_backward_workspace_bytes(a.rows, a.in_features, a.out_features);
        if (size > 0) {
          work = at::empty({size}, options.dtype(at::kByte));
          a.workspace = work.data_ptr();
          a.workspace_bytes = size;
        }
        check_call("rfm_linear_backward", rfm_linear_backward(&a, current_stream(dy.device())));
      }
    }
    return once(std::move(result), "linear");
  }
};

// Under autocast the operands take its type, as torch's own linear does.
Tensor lowered(const Tensor& t, at::ScalarType type) {
  return t.defined() && t.is_floating_point() && t.scalar_type() != at::kDouble && t.scalar_type() != type
             ? t.to(type)
             : t;
}

}  // namespace

Tensor linear(const Tensor& x_in, const Tensor& weight_in, const MaybeTensor& maybe_bias, int64_t activation,
              const MaybeTensor& maybe_residual) {
  refuse_traced("linear");
  Tensor x = x_in, weight = weight_in, bias = or_undefined(maybe_bias), residual = or_undefined(maybe_residual);
  refuse_tangents("linear", {&x, &weight, &bias, &residual});
  RFM_REQUIRE(x.is_cuda(), "x must be a CUDA tensor (linear has no CPU path)");
  RFM_REQUIRE(activation >= RFM_ACT_NONE && activation <= RFM_ACT_GELU, "unknown activation ", activation);
  RFM_REQUIRE(weight.dim() == 2 && weight.device() == x.device(), "weight must be a matrix on x's device");
  const int64_t in = weight.size(1), out = weight.size(0);
  RFM_REQUIRE(in >= 1 && out >= 1 && in <= (1 << 30) && out <= (1 << 30),
              "weight must have at least one row and one column");
  RFM_REQUIRE(x.dim() >= 1 && x.size(-1) == in, "x must end in a dimension of ", in, " like weight's rows, got ",
              x.sizes());
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {
    const at::ScalarType type = at::autocast::get_autocast_dtype(at::kCUDA);
    x = lowered(x, type);
    weight = lowered(weight, type);
    residual = lowered(residual, type);
    if (bias.defined() && bias.scalar_type() != at::kFloat) bias = lowered(bias, type);
  }
  RFM_REQUIRE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
              "x must be bfloat16 or float16 (the tensor cores' types), got ", x.scalar_type());
  RFM_REQUIRE(weight.scalar_type() == x.scalar_type(), "weight must have x's type, got ", weight.scalar_type());
  if (bias.defined()) {
    RFM_REQUIRE(bias.device() == x.device() && bias.dim() == 1 && bias.size(0) == out, "bias must have shape [", out,
                "] on x's device");
    RFM_REQUIRE(bias.scalar_type() == x.scalar_type() || bias.scalar_type() == at::kFloat,
                "bias must be float32 or of x's type, got ", bias.scalar_type());
    if (!bias.is_contiguous()) bias = bias.contiguous();
  }
  if (residual.defined()) {
    RFM_REQUIRE(residual.device() == x.device() && residual.scalar_type() == x.scalar_type(),
                "residual must have x's type and device");
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = out;
    RFM_REQUIRE(residual.sizes() == at::IntArrayRef(shape), "residual must have the output's shape ",
                at::IntArrayRef(shape), ", got ", residual.sizes());
  }
  const c10::cuda::CUDAGuard guard(x.device());
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual))) {
    return Linear::apply(x, weight, maybe(bias), activation, maybe(residual));
  }
  return forward_rows(x, weight, bias, activation, residual, false).out;
}

}  // namespace rfm_host
