// layer_norm: checks, allocation and autograd around rfm_layer_norm_*.
#include "host_common.h"

namespace rfm_host {
namespace {

struct Outputs {
  Tensor out, stats;
};

int param_code(const Tensor& x, const Tensor& weight, const Tensor& bias) {
  const Tensor& p = weight.defined() ? weight : bias;
  return dtype_code(p.defined() ? p.scalar_type() : x.scalar_type());
}

Outputs forward_rows(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, bool stats) {
  Outputs o;
  const Tensor rows = rows_of(x);
  const int64_t n = rows.size(0), dim = rows.size(1);
  o.out = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  if (stats) o.stats = at::empty({2, n}, x.options().dtype(at::kFloat));
  if (n > 0) {
    float* mean = stats ? o.stats.data_ptr<float>() : nullptr;
    check_call("rfm_layer_norm_forward",
               rfm_layer_norm_forward(rows.data_ptr(), row_stride(rows), data_or_null(weight), data_or_null(bias),
                                      o.out.data_ptr(), mean, stats ? mean + n : nullptr, n, static_cast<int>(dim),
                                      static_cast<float>(eps), dtype_code(x.scalar_type()),
                                      param_code(x, weight, bias), current_stream(x.device())));
  }
  return o;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& maybe_weight,
                        const MaybeTensor& maybe_bias, double eps) {
    const Tensor weight = or_undefined(maybe_weight), bias = or_undefined(maybe_bias);
    at::AutoDispatchBelowADInplaceOrView guard;
    Outputs o = forward_rows(x, weight, bias, eps, true);
    // x itself, not a view made here: only it shares the version that an in-place change advances
    ctx->save_for_backward({x, weight, o.stats});
    ctx->saved_data["param"] = static_cast<int64_t>(param_code(x, weight, bias));
    // places among the tensors given (-1: not given), which number the gradients asked for
    ctx->saved_data["weight"] = static_cast<int64_t>(weight.defined() ? 1 : -1);
    ctx->saved_data["bias"] = static_cast<int64_t>(bias.defined() ? (weight.defined() ? 2 : 1) : -1);
    return o.out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    refuse_tangents("layer_norm's gradient", {&grads[0]});
    const Tensor& x = saved[0];
    // saved-tensor hooks may have given everything other strides
    const Tensor weight = saved[1].defined() ? saved[1].contiguous() : Tensor(), stats = saved[2].contiguous();
    const c10::cuda::CUDAGuard guard(x.device());
    variable_list result(4);
    {
      at::AutoGradMode off(false);
      const Tensor rows = rows_of(x);
      const int64_t n = rows.size(0), dim = rows.size(1);
      const int64_t param = ctx->saved_data["param"].toInt();
      const auto kind = param == RFM_DTYPE_F32 ? at::kFloat : param == RFM_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
      const Tensor g = rows_of(grads[0].scalar_type() == rows.scalar_type() ? grads[0]
                                                                            : grads[0].to(rows.scalar_type()));
      if (ctx->needs_input_grad(0)) {
        result[0] = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
      }
      const int64_t at_w = ctx->saved_data["weight"].toInt(), at_b = ctx->saved_data["bias"].toInt();
      if (at_w > 0 && ctx->needs_input_grad(at_w)) result[1] = at::empty({dim}, rows.options().dtype(kind));
      if (at_b > 0 && ctx->needs_input_grad(at_b)) result[2] = at::empty({dim}, rows.options().dtype(kind));
      int64_t size = 0;
      Tensor work;
      if (result[1].defined() || result[2].defined()) {
        size = rfm_layer_norm_workspace_bytes(n, static_cast<int>(dim));
        if (size > 0) work = at::empty({size}, rows.options().dtype(at::kByte));
      }
      const float* mean = stats.data_ptr<float>();
      check_call("rfm_layer_norm_backward",
                 rfm_layer_norm_backward(rows.data_ptr(), row_stride(rows), data_or_null(weight), mean, mean + n,
                                         g.data_ptr(), row_stride(g), data_or_null(result[0]),
                                         data_or_null(result[1]), data_or_null(result[2]), n, static_cast<int>(dim),
                                         dtype_code(rows.scalar_type()), static_cast<int>(param), data_or_null(work),
                                         size, current_stream(rows.device())));
    }
    return once(std::move(result), "layer_norm");
  }
};

}  // namespace

Tensor layer_norm(const Tensor& x, const MaybeTensor& maybe_weight, const MaybeTensor& maybe_bias, double eps) {
  refuse_traced("layer_norm");
  Tensor weight = or_undefined(maybe_weight), bias = or_undefined(maybe_bias);
  refuse_tangents("layer_norm", {&x, &weight, &bias});
  RFM_REQUIRE(x.is_cuda(), "x must be a CUDA tensor (layer_norm has no CPU path)");
  RFM_REQUIRE(dtype_code(x.scalar_type()) >= 0, "x must be float32, bfloat16 or float16, got ", x.scalar_type());
  RFM_REQUIRE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= (1 << 30),
              "x needs a last dimension of at least one element");
  RFM_REQUIRE(eps >= 0.0, "eps must not be negative, got ", eps);
  for (const Tensor* p : {&weight, &bias}) {
    if (!p->defined()) continue;
    const char* name = p == &weight ? "weight" : "bias";
    RFM_REQUIRE(p->device() == x.device() && p->dim() == 1 && p->size(0) == x.size(-1), name, " must have shape [",
                x.size(-1), "] on x's device");
    RFM_REQUIRE(p->scalar_type() == x.scalar_type() || p->scalar_type() == at::kFloat, name,
                " must be float32 or of x's type, got ", p->scalar_type());
  }
  RFM_REQUIRE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
              "weight and bias must have one type");
  if (weight.defined() && !weight.is_contiguous()) weight = weight.contiguous();
  if (bias.defined() && !bias.is_contiguous()) bias = bias.contiguous();
  const c10::cuda::CUDAGuard guard(x.device());
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias))) {
    return LayerNorm::apply(x, maybe(weight), maybe(bias), eps);
  }
  return forward_rows(x, weight, bias, eps, false).out;
}

}  // namespace rfm_host
